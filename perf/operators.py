"""Measured cases of the language-model operators around the scans: the residual
RMSNorm with an int8 output, the int8 linear layer, and the gated linear
recurrence with its backward pass and single-token step.

``run`` computes a case either with the package's operators (``own`` true) or
with elementary torch operations in 32 bits (``own`` false); ``exact`` gives the
same outputs from the definitions in 64 bits.

Definitions
    add_rmsnorm        s = x + residual in the residual's type, y = w s / sqrt(mean(s^2) + eps)
    ..._int8           scale = max|y| / 127 per row, q = rint(y / scale)
    int8_linear        y[m, n] = scale[m] wscale[n] sum_k q[m, k] wq[n, k] + bias[n]
    gated recurrence   g_t = (1 - lower) sigmoid(-forget_t)
                       h_t = (1 - g_t) h_{t-1} + g_t x_t      (h_{t-1} = 0 where reset_t)
                       y_t = h_t silu(z_t)
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5


def listed():
    return [
        # one decode step of eight sequences: the latency of the norm in front of a projection
        dict(name="norm_int8_decode", op="norm_int8", rows=8, features=2560, dtype="bf16", residual=True),
        # a prompt batch of two 8192-token sequences at the Mamba-2 layer's width
        dict(name="norm_int8_prefill", op="norm_int8", rows=16384, features=2560, dtype="bf16", residual=True),
        # an odd width whose rows have no 16-byte alignment, first layer (no residual yet)
        dict(name="norm_int8_odd", op="norm_int8", rows=1031, features=2051, dtype="f16", residual=False),
        # the training step of the pre-norm at the layer's 8 x 8192 tokens, residual stream in 32 bits
        dict(name="norm_train", op="norm_train", rows=65536, features=2560, dtype="bf16", residual=True),
        # the in-projection of one token: reading the weights once is all there is
        dict(name="linear_token", op="linear", m=1, k=2560, n=12368, dtype="bf16", bias=False, dynamic=False),
        # the out-projection of a decode batch, activations quantised in the same pass
        dict(name="linear_batch", op="linear", m=100, k=5120, n=2560, dtype="bf16", bias=True, dynamic=True),
        # the in-projection of a ragged prompt of 1531 tokens, half precision out
        dict(name="linear_ragged", op="linear", m=1531, k=2560, n=12368, dtype="f16", bias=True, dynamic=False),
        # the in-projection of 8 x 8192 prompt tokens
        dict(name="linear_prefill", op="linear", m=65536, k=2560, n=12368, dtype="bf16", bias=False, dynamic=False),
        # one decode step of 128 sequences
        dict(name="recurrence_step", op="step", batch=128, dim=5120, dtype="bf16", gate=True),
        # one 4096-token prompt: few rows, so the sequence has to be cut
        dict(name="recurrence_prompt", op="scan", batch=1, length=4096, dim=5120, dtype="bf16", gate=True, packed=False),
        # training on three packed rows of odd length, odd width and 32-bit storage
        dict(name="recurrence_packed", op="scan_train", batch=3, length=5003, dim=1283, dtype="f32", gate=False,
             packed=True),
        # training at the selective scan's headline shape
        dict(name="recurrence_train", op="scan_train", batch=16, length=4096, dim=5120, dtype="bf16", gate=True,
             packed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_int8", "norm_train", "linear", "linear", "step", "scan", "scan_train"])
    if op.startswith("norm"):
        features = _log(rng, 256, 8192)
        if rng.random() < 0.7:
            features = max(256, features // 64 * 64)
        rows = min(_log(rng, 1, 65536), 65536 * 2560 // features)
        dtype = "bf16" if op == "norm_train" else rng.choice(["bf16", "f16"])
        return dict(op=op, rows=rows, features=features, dtype=dtype,
                    residual=op == "norm_train" or rng.random() < 0.7)
    if op == "linear":
        k, n = _log(rng, 256, 8192), _log(rng, 256, 16384)
        if rng.random() < 0.75:
            k, n = max(256, k // 16 * 16), max(256, n // 16 * 16)
        m = min(_log(rng, 1, 65536), 65536 * 2560 * 12368 // (k * n))
        return dict(op=op, m=m, k=k, n=n, dtype=rng.choice(["bf16", "f16"]), bias=rng.random() < 0.5,
                    dynamic=rng.random() < 0.5)
    dim = _log(rng, 96, 8192)
    if rng.random() < 0.7:
        dim = max(96, dim // 32 * 32)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "step":
        return dict(op=op, batch=_log(rng, 1, 1024), dim=dim, dtype=dtype, gate=rng.random() < 0.7)
    top = 16 * 4096 * 5120 // (2 if dtype == "f32" else 1)
    batch = _log(rng, 1, 16)
    length = min(_log(rng, 1, 65536), top // (dim * batch))
    return dict(op=op, batch=batch, length=length, dim=dim, dtype=dtype, gate=rng.random() < 0.6,
                packed=rng.random() < 0.4)


# ------------------------------------------------------------------ inputs --
def _rows_int8(t):
    """Weights and activations as a checkpoint or an earlier layer leaves them: int8 rows and their scales."""
    scale = t.abs().amax(dim=1) / 127.0
    return torch.round(t / scale[:, None]).clamp_(-127, 127).to(torch.int8), scale


def _activations(g, rows, features, dtype):
    """Unit normal with a few channels of large values, as residual streams have them."""
    x = torch.randn(rows, features, device="cuda", generator=g, dtype=torch.float32 if dtype == "f32" else _DT[dtype])
    x[:, :: max(1, features // 5)] *= 8
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    dt = _DT[case["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    s = dict(case=case)
    if op.startswith("norm"):
        rows, features = case["rows"], case["features"]
        train = op == "norm_train"
        s["x"] = _activations(g, rows, features, case["dtype"])
        s["residual"] = randn(rows, features, dtype=torch.float32 if train else dt) if case["residual"] else None
        s["weight"] = 1 + 0.1 * randn(features)
        if train:
            s["dy"] = randn(rows, features, dtype=dt)
            s["ds"] = randn(rows, features)
            for k in ("x", "residual", "weight"):
                s[k].requires_grad_(True)
    elif op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        if case["dynamic"]:
            s["x"] = _activations(g, m, k, case["dtype"])
        else:
            s["q"], s["scale"] = _rows_int8(randn(m, k, dtype=torch.float16).float())
        s["wq"], s["wscale"] = _rows_int8(randn(n, k) / math.sqrt(k))
        s["bias"] = 0.1 * randn(n) if case["bias"] else None
    else:
        batch, dim = case["batch"], case["dim"]
        shape = (batch, dim) if op == "step" else (batch, case["length"], dim)
        s["x"] = randn(*shape, dtype=dt)
        s["forget"] = randn(*shape, dtype=dt).mul_(1.5).add_(2.0)     # gates that mostly keep their state
        s["z"] = randn(*shape, dtype=dt) if case["gate"] else None
        s["lower"] = torch.rand(dim, device="cuda", generator=g) * 0.9
        s["state"] = randn(batch, dim)
        if op != "step":
            s["reset"] = (torch.rand(batch, case["length"], device="cuda", generator=g) < 1 / 700) \
                if case["packed"] else None
        if op == "scan_train":
            s["dy"] = randn(*shape, dtype=dt)
            s["dstate"] = randn(batch, dim)
            for k in ("x", "forget", "z", "lower", "state"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------- the operators --
def _values(q, scale, dtype):
    """What int8 rows stand for, in the activations' type."""
    return torch.mul(q, scale[..., None], out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _run_own(s):
    from metal_kernelops_b200 import cv
    c = s["case"]
    op, dt = c["op"], _DT[c["dtype"]]
    if op == "norm_int8":
        q, scale, stream = cv.add_rmsnorm_int8(s["x"], s["weight"], s["residual"], eps=EPS)
        return dict(y=_values(q, scale, dt), scale=scale, stream=stream)
    if op == "norm_train":
        y, stream = cv.add_rmsnorm(s["x"], s["weight"], s["residual"], eps=EPS)
        dx, dres, dw = torch.autograd.grad((y, stream), (s["x"], s["residual"], s["weight"]), (s["dy"], s["ds"]))
        return dict(y=y.detach(), stream=stream.detach(), dx=dx, dres=dres, dweight=dw)
    if op == "linear":
        q, scale = cv.quantize_int8(s["x"]) if c["dynamic"] else (s["q"], s["scale"])
        return cv.int8_linear(q, scale, s["wq"], s["wscale"], s["bias"], out_dtype=dt)
    if op == "step":
        y = cv.gated_linear_recurrence_update(s["state"], s["x"], s["forget"], s["z"], lower_bound=s["lower"])
        return dict(y=y, state=s["state"])
    if op == "scan":
        with torch.no_grad():
            y, final = cv.gated_linear_recurrence(s["x"], s["forget"], s["z"], lower_bound=s["lower"],
                                                  initial_state=s["state"], reset=s["reset"])
        return dict(y=y, final=final)
    y, final = cv.gated_linear_recurrence(s["x"], s["forget"], s["z"], lower_bound=s["lower"],
                                          initial_state=s["state"], reset=s["reset"])
    names = [k for k in ("x", "forget", "z", "lower", "state") if s[k] is not None]
    grads = torch.autograd.grad((y, final), [s[k] for k in names], (s["dy"], s["dstate"]))
    return dict(y=y.detach(), final=final.detach(), **{"d" + k: v for k, v in zip(names, grads)})


# ------------------------------------------------------------ plain forms --
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, doubling the span a step at a time; overwrites a and b."""
    span, length = 1, a.shape[1]
    while span < length:
        b[:, span:] += a[:, span:] * b[:, :-span]
        a[:, span:] = a[:, span:] * a[:, :-span]
        span *= 2
    return b


def _plain_norm(s):
    c = s["case"]
    dt = _DT[c["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    stream = x if s["residual"] is None else x + s["residual"].float()
    kept = stream.to(s["x"].dtype if s["residual"] is None else s["residual"].dtype)
    h = kept.float()
    rstd = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
    xh = h * rstd
    y = xh * w
    if c["op"] == "norm_int8":
        scale = y.abs().amax(dim=1) / 127.0
        q = torch.round(y / scale[:, None]).to(torch.int8)
        return dict(y=_values(q, scale, dt), scale=scale, stream=kept)
    dy = s["dy"].float()
    dxh = dy * w
    d = rstd * (dxh - xh * (dxh * xh).mean(dim=1, keepdim=True)) + s["ds"]
    return dict(y=y.to(dt), stream=kept, dx=d.to(dt), dres=d, dweight=(dy * xh).sum(dim=0))


def _plain_linear(s):
    c = s["case"]
    if c["dynamic"]:
        x = s["x"].float()
        scale = x.abs().amax(dim=1) / 127.0
        q = torch.round(x / scale[:, None])
    else:
        q, scale = s["q"].float(), s["scale"]
    y = torch.matmul(q, s["wq"].float().t())
    y = y * scale[:, None] * s["wscale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(_DT[c["dtype"]])


def _plain_scan(s):
    c = s["case"]
    dt = _DT[c["dtype"]]
    x, forget, span = s["x"].float(), s["forget"].float(), 1 - s["lower"]
    keep_in = torch.sigmoid(-forget)
    g = span * keep_in
    if c["op"] == "step":
        h = s["state"] + g * (x - s["state"])
        y = h if s["z"] is None else h * (s["z"].float() * torch.sigmoid(s["z"].float()))
        return dict(y=y.to(dt), state=s["state"].copy_(h))      # in place, as a decode loop keeps it
    a = 1 - g
    if s["reset"] is not None:
        a = a.masked_fill(s["reset"][..., None], 0.0)
    b = g * x
    b[:, 0] += a[:, 0] * s["state"]
    h = _scan(a.clone(), b)
    if s["z"] is None:
        sg = None
        y = h.to(dt)
    else:
        z = s["z"].float()
        sg = torch.sigmoid(z)
        y = (h * (z * sg)).to(dt)
    out = dict(y=y, final=h[:, -1].clone())
    if c["op"] == "scan":
        return out
    dy = s["dy"].float()
    if sg is not None:
        out["dz"] = (dy * h * (sg * (1 + z * (1 - sg)))).to(dt)
        dy = dy * (z * sg)
        del z, sg
    before = torch.cat([s["state"][:, None], h[:, :-1]], dim=1)
    if s["reset"] is not None:
        before = before.masked_fill(s["reset"][..., None], 0.0)
    first = a[:, 0].clone()
    # dh_t = dy_t + a_{t+1} dh_{t+1}: the same scan over the reversed sequence
    back = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], dim=1).flip(1)
    del a, h, b
    dh = dy.flip(1)
    dh[:, 0] += s["dstate"]
    back[:, 0] = 0.0
    dh = _scan(back, dh).flip(1)
    out["dx"] = (g * dh).to(dt)
    dg = dh * (x - before)
    out["dforget"] = (-dg * g * torch.sigmoid(forget)).to(dt)
    out["dlower"] = -(dg * keep_in).sum(dim=(0, 1))
    out["dstate"] = first * dh[:, 0]
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        if op.startswith("norm"):
            return _plain_norm(state)
        return _plain_linear(state) if op == "linear" else _plain_scan(state)


# --------------------------------------------------------------- the work --
def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op.startswith("norm"):
        n = case["rows"] * case["features"]
        if op == "norm_int8":
            per = (3 * e if case["residual"] else e) + 1     # x, residual -> stream, int8; without a residual x is the stream
            return {"bytes": n * per + 4 * (case["rows"] + case["features"]), "flops": 8 * n}
        # forward x, residual -> stream, y; backward stream, dy, dstream -> dx, dresidual
        return {"bytes": n * ((e + 4 + 4 + e) + (4 + e + 4 + e + 4)) + 8 * case["features"], "flops": 20 * n}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        inp = m * k * (e if case["dynamic"] else 1) + (0 if case["dynamic"] else 4 * m)
        return {"bytes": inp + n * k + 4 * n + (4 * n if case["bias"] else 0) + m * n * e, "flops": 2 * m * k * n}
    tensors = 3 if case["gate"] else 2
    if op == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (e * (tensors + 1) + 8) + 4 * case["dim"], "flops": 20 * n}
    n = case["batch"] * case["length"] * case["dim"]
    fixed = 8 * case["batch"] * case["dim"] + 4 * case["dim"] + (case["batch"] * case["length"] if case["packed"] else 0)
    if op == "scan":
        return {"bytes": n * e * (tensors + 1) + fixed, "flops": 20 * n}
    return {"bytes": n * e * ((tensors + 1) + (2 * tensors + 1)) + 3 * fixed, "flops": 60 * n}


# ------------------------------------------------------- 64-bit definitions --
def _exact_norm(s):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    if s["residual"] is None:
        h = x
    else:
        h = (x + s["residual"].detach().double()).to(s["residual"].dtype).double()
    ms = torch.einsum("rf,rf->r", h, h) / h.shape[1] + EPS
    n = h / torch.sqrt(ms)[:, None]
    y = n * w[None]
    if s["case"]["op"] == "norm_int8":
        scale = y.abs().max(dim=1).values / 127
        return dict(y=torch.round(y / scale[:, None]) * scale[:, None], scale=scale, stream=h)
    up = s["dy"].double()
    inner = torch.einsum("rf,rf,f->r", up, n, w) / h.shape[1]
    d = (up * w[None] - n * inner[:, None]) / torch.sqrt(ms)[:, None] + s["ds"].double()
    return dict(y=y, stream=h, dx=d, dres=d, dweight=torch.einsum("rf,rf->f", up, n))


def _exact_linear(s):
    if s["case"]["dynamic"]:
        x = s["x"].double()
        scale = x.abs().max(dim=1).values / 127
        q = torch.round(x / scale[:, None])
    else:
        q, scale = s["q"].double(), s["scale"].double()
    y = torch.nn.functional.linear(q * scale[:, None], s["wq"].double() * s["wscale"].double()[:, None])
    return y if s["bias"] is None else y.add_(s["bias"].double())


def _exact_scan(s):
    c = s["case"]
    one = c["op"] == "step"
    x, forget, z = (None if s[k] is None else s[k].detach().double() for k in ("x", "forget", "z"))
    if one:
        x, forget, z = (None if t is None else t[:, None] for t in (x, forget, z))
    lower = s["lower"].detach().double()
    state = s["state"].detach().double()
    reset = None if one else s["reset"]
    length = x.shape[1]
    f = lower + (1 - lower) / (1 + torch.exp(-forget))
    g = (1 - lower) / (1 + torch.exp(forget))
    past = torch.empty_like(x)          # the state that enters each step, zero after a reset
    hs = torch.empty_like(x)
    h = state
    for t in range(length):
        if reset is not None:
            h = torch.where(reset[:, t, None], torch.zeros_like(h), h)
        past[:, t] = h
        h = torch.addcmul(f[:, t] * h, g[:, t], x[:, t])
        hs[:, t] = h
    gate = None if z is None else z / (1 + torch.exp(-z))
    y = hs if gate is None else hs * gate
    if one:
        return dict(y=y[:, 0], state=h)
    out = dict(y=y, final=h)
    if c["op"] == "scan":
        return out
    up = s["dy"].double()
    if gate is not None:
        sz = 1 / (1 + torch.exp(-z))
        out["dz"] = up * hs * (sz + gate * (1 - sz))
        up = up * gate
        del sz, gate
    del hs, y
    dh = torch.empty_like(x)
    d = s["dstate"].double()
    for t in range(length - 1, -1, -1):
        d = d + up[:, t]
        dh[:, t] = d
        d = d * f[:, t]
        if reset is not None:
            d = torch.where(reset[:, t, None], torch.zeros_like(d), d)
    df = dh.mul(past - x)               # h = f past + (1 - f) x
    out["dx"] = dh * g
    sig = 1 / (1 + torch.exp(-forget))
    out["dforget"] = df * ((1 - lower) * sig * (1 - sig))
    out["dlower"] = (df * (1 - sig)).sum(dim=(0, 1))
    out["dstate"] = d
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("scan", "scan_train") and case["length"] > 100000:
        return None
    with torch.no_grad():
        if case["op"].startswith("norm"):
            return _exact_norm(s)
        return _exact_linear(s) if case["op"] == "linear" else _exact_scan(s)
