"""The language-model operators under tracers, dispatch modes, transforms and the compiler.

Whatever records or rewrites a program has to see each call as its registered operator: a
recorded graph that holds an allocation in the place of the call would return memory that
nothing wrote.  All comparisons are bit for bit: the same kernels run on the same values.
"""

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _cv():
    from metal_kernelops_b200 import cv
    return cv


def _ops(device="cuda"):
    """name -> (registered operator, function of tensors, its tensors)."""
    cv = _cv()
    g = torch.Generator().manual_seed(1)

    def r(*shape, dtype=F32):
        return torch.randn(*shape, generator=g).to(device, dtype)

    x, w, res = r(6, 64, dtype=BF16), 1 + 0.1 * r(64), r(6, 64)
    q = torch.randint(-127, 128, (6, 64), generator=g, dtype=torch.int8).to(device)
    wq = torch.randint(-127, 128, (24, 64), generator=g, dtype=torch.int8).to(device)
    qs, ws = torch.rand(6, generator=g).to(device), torch.rand(24, generator=g).to(device)
    sx, sf, sz = r(2, 70, 64, dtype=BF16), r(2, 70, 64, dtype=BF16), r(2, 70, 64, dtype=BF16)

    def step(state, x, f, z):
        state = state.clone()
        return cv.gated_linear_recurrence_update(state, x, f, z), state

    return {
        "add_rmsnorm": ("add_rmsnorm_fwd", lambda x, w, res: cv.add_rmsnorm(x, w, res), (x, w, res)),
        "add_rmsnorm_int8": ("add_rmsnorm_int8", lambda x, w, res: cv.add_rmsnorm_int8(x, w, res), (x, w, res)),
        "quantize_int8": ("quantize_int8", cv.quantize_int8, (x,)),
        "int8_linear": ("int8_linear", lambda q, qs, wq, ws: cv.int8_linear(q, qs, wq, ws), (q, qs, wq, ws)),
        "recurrence": ("gated_recurrence_fwd", lambda x, f, z: cv.gated_linear_recurrence(x, f, z), (sx, sf, sz)),
        "update": ("gated_recurrence_update", step, (r(2, 64), sx[:, 0], sf[:, 0], sz[:, 0])),
    }


NAMES = ["add_rmsnorm", "add_rmsnorm_int8", "quantize_int8", "int8_linear", "recurrence", "update"]


def _flat(out):
    return [out] if isinstance(out, torch.Tensor) else list(out)


def _other(ts):
    """Other values of the same shapes."""
    g = torch.Generator(device="cuda").manual_seed(2)
    return [torch.randint(-127, 128, t.shape, device="cuda", dtype=torch.int8, generator=g) if t.dtype == torch.int8
            else (torch.randn(t.shape, device="cuda", generator=g).abs() + 0.1).to(t.dtype) for t in ts]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@torch.no_grad()
def test_make_fx_records_the_operator(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    op, fn, ts = _ops()[name]
    graph = make_fx(fn)(*ts)
    assert any(op in str(n.target) for n in graph.graph.nodes)
    new = _other(ts)
    assert all(torch.equal(a, b) for a, b in zip(_flat(graph(*new)), _flat(fn(*new))))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.filterwarnings("ignore")
@torch.no_grad()
def test_jit_trace_records_the_operator(name):
    op, fn, ts = _ops()[name]
    traced = torch.jit.trace(lambda *a: tuple(_flat(fn(*a))), tuple(ts), check_trace=False)
    assert op in str(traced.graph)
    new = _other(ts)
    assert all(torch.equal(a, b) for a, b in zip(traced(*new), _flat(fn(*new))))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@torch.no_grad()
def test_dispatch_modes_see_the_operator(name):
    from torch.utils._python_dispatch import TorchDispatchMode
    op, fn, ts = _ops()[name]
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Log():
        out = fn(*ts)
    assert any(op in s for s in seen)
    assert all(torch.equal(a, b) for a, b in zip(_flat(out), _flat(fn(*ts))))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["add_rmsnorm", "add_rmsnorm_int8", "quantize_int8", "int8_linear", "recurrence"])
@pytest.mark.filterwarnings("ignore")
@torch.no_grad()
def test_vmap(name):
    _, fn, ts = _ops()[name]
    many = [_other(ts), list(ts), _other(ts)]
    got = torch.vmap(fn)(*(torch.stack(t) for t in zip(*many)))
    for i, one in enumerate(many):
        assert all(torch.equal(a[i], b) for a, b in zip(_flat(got), _flat(fn(*one))))


@pytest.mark.gpu
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_training(dynamic):
    """torch.compile of a layer with its gradients, at two lengths."""
    cv = _cv()

    def layer(x, w, res, forget, z):
        y, stream = cv.add_rmsnorm(x, w, res)
        y, final = cv.gated_linear_recurrence(y, forget, z)
        return y.float().sum() + (stream * stream).sum() + final.sum()

    compiled = torch.compile(layer, fullgraph=True, backend="aot_eager", dynamic=dynamic)
    g = torch.Generator(device="cuda").manual_seed(1)
    for length in (5, 70):
        x, forget, z = (torch.randn(2, length, 64, device="cuda", generator=g).to(BF16).requires_grad_(True)
                        for _ in range(3))
        res = torch.randn(2, length, 64, device="cuda", generator=g).requires_grad_(True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        leaves = (x, w, res, forget, z)
        a, b = (torch.autograd.grad(fn(*leaves), leaves) for fn in (compiled, layer))
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dynamic", [False, True])
@torch.no_grad()
def test_compiled_serving(dynamic):
    """torch.compile of a decode step: the state is updated in place."""
    cv = _cv()

    def token(x, w, res, wq, ws, forget, state):
        q, scale, stream = cv.add_rmsnorm_int8(x, w, res)
        h = cv.int8_linear(q, scale, wq, ws)
        y = cv.gated_linear_recurrence_update(state, h, forget)
        return (*cv.quantize_int8(y), stream)

    compiled = torch.compile(token, fullgraph=True, backend="aot_eager", dynamic=dynamic)
    g = torch.Generator(device="cuda").manual_seed(1)
    wq, ws = cv.quantize_int8(torch.randn(32, 64, device="cuda", generator=g))
    for batch in (5, 9):
        x = torch.randn(batch, 64, device="cuda", generator=g).to(BF16)
        res, w = torch.randn(batch, 64, device="cuda", generator=g), torch.ones(64, device="cuda")
        forget = torch.randn(batch, 32, device="cuda", generator=g).to(BF16)
        s1 = torch.randn(batch, 32, device="cuda", generator=g)
        s2 = s1.clone()
        a, b = compiled(x, w, res, wq, ws, forget, s1), token(x, w, res, wq, ws, forget, s2)
        assert all(torch.equal(u, v) for u, v in zip(a, b)) and torch.equal(s1, s2)


@pytest.mark.gpu
def test_registered_operators_pass_opcheck():
    ops = torch.ops.b200ssm
    g = torch.Generator(device="cuda").manual_seed(1)

    def r(*shape, grad=False):
        return torch.randn(*shape, device="cuda", generator=g).requires_grad_(grad)

    q, wq = torch.ones(5, 64, dtype=torch.int8, device="cuda"), torch.ones(8, 64, dtype=torch.int8, device="cuda")
    reset = torch.zeros(2, 5, dtype=torch.bool, device="cuda")
    for op, args in (
            (ops.add_rmsnorm_fwd, (r(5, 64, grad=True), r(64, grad=True), r(5, 64, grad=True), 1e-5, True)),
            (ops.add_rmsnorm_fwd, (r(5, 64, grad=True), r(64, grad=True), None, 1e-5, True)),
            (ops.add_rmsnorm_int8, (r(5, 64), r(64), r(5, 64), 1e-5)),
            (ops.int8_linear, (q, r(5), wq, r(8), None, F16)),
            (ops.gated_recurrence_fwd, (*(r(2, 5, 64, grad=True) for _ in range(3)), torch.rand(64, device="cuda"),
                                        r(2, 64, grad=True), reset, True)),
            (ops.gated_recurrence_update, (r(2, 64), r(2, 64), r(2, 64), r(2, 64), r(64)))):
        torch.library.opcheck(op.default, args)


# --------------------------------------------------------------- without a GPU --
def test_direct_calls_step_aside_for_whatever_watches(monkeypatch):
    """The choice itself, on CPU tensors that stand for tensors of the current device."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    from metal_kernelops_b200 import _native as nat
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    x = torch.ones(2)
    assert nat.direct(x, None, torch.nn.Parameter(x))
    seen = []

    def note(t):
        seen.append(nat.direct(t))
        return t + 1

    make_fx(note)(x)
    torch.jit.trace(note, (x,), check_trace=False)
    torch.vmap(note)(x)
    torch.func.grad(lambda t: note(t).sum())(x)

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Mode():
        note(x)
    with FakeTensorMode():
        seen.append(nat.direct(x))
    assert seen and not any(seen)
    assert nat.direct(x)
