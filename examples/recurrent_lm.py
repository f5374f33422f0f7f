"""A small recurrent language model on the package's operators: trained in bfloat16,
then served in 8-bit integers.

    python examples/recurrent_lm.py [--layers 4] [--width 512] [--steps 60]

A layer is ``stream = stream + out(recurrence(in(norm(stream))))``:

* training: ``add_rmsnorm`` (the residual's addition and the norm in one pass, the
  stream in float32), the projections in bfloat16, ``gated_linear_recurrence`` with
  its backward pass over packed sequences;
* serving: ``add_rmsnorm_int8`` hands int8 rows to ``int8_linear``, the recurrence runs
  the prompt and keeps its state, ``quantize_int8`` prepares the out-projection's
  input, and ``gated_linear_recurrence_update`` takes one token per sequence; the
  decode step is captured in a CUDA graph.

The data are synthetic: sequences that repeat a random motif, so that a model with
memory beats one without.
"""

from __future__ import annotations

import argparse
import pathlib
import sys
import time

import torch
import torch.nn.functional as F

ROOT = pathlib.Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from metal_kernelops_b200 import check_errors, cv  # noqa: E402


class Layer(torch.nn.Module):
    def __init__(self, width, inner, depth):
        super().__init__()
        self.inner = inner
        self.norm = torch.nn.Parameter(torch.ones(width))
        self.in_proj = torch.nn.Linear(width, 3 * inner)            # x, forget gate, output gate
        self.out_proj = torch.nn.Linear(inner, width)
        self.lower = torch.nn.Parameter(torch.full((inner,), depth))  # deeper layers remember longer
        with torch.no_grad():
            self.in_proj.bias[inner:2 * inner].uniform_(0.0, 4.0)

    def lower_bound(self):
        return self.lower.clamp(0.0, 0.99)

    def forward(self, h, stream, reset):
        """h: the previous layer's output, joined to the stream here."""
        y, stream = cv.add_rmsnorm(h, self.norm, stream)
        x, forget, z = F.linear(y, self.in_proj.weight.to(y.dtype), self.in_proj.bias.to(y.dtype)).split(self.inner, -1)
        y, _ = cv.gated_linear_recurrence(x, forget, z, lower_bound=self.lower_bound(), reset=reset)
        return F.linear(y, self.out_proj.weight.to(y.dtype), self.out_proj.bias.to(y.dtype)), stream


class Model(torch.nn.Module):
    def __init__(self, vocab=64, width=512, inner=768, layers=4):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width)
        self.layers = torch.nn.ModuleList(Layer(width, inner, 0.9 * i / max(1, layers - 1)) for i in range(layers))
        self.norm = torch.nn.Parameter(torch.ones(width))
        self.head = torch.nn.Linear(width, vocab, bias=False)

    def forward(self, tokens, reset=None):
        """Logits (batch, length, vocab) in float32."""
        stream = self.embed(tokens).float()
        h = torch.zeros(stream.shape, dtype=torch.bfloat16, device=stream.device)
        for layer in self.layers:
            h, stream = layer(h, stream, reset)
        y, _ = cv.add_rmsnorm(h, self.norm, stream)
        return F.linear(y, self.head.weight.to(y.dtype)).float()


class Served:
    """The model's weights in int8, one scale per output feature."""

    @torch.no_grad()
    def __init__(self, model):
        def quantised(linear):
            return (*cv.quantize_int8(linear.weight), None if linear.bias is None else linear.bias.clone())

        self.embed = model.embed.weight.float().clone()
        self.layers = [dict(norm=m.norm.clone(), inner=m.inner, lower=m.lower_bound(),
                            proj_in=quantised(m.in_proj), proj_out=quantised(m.out_proj)) for m in model.layers]
        self.norm, self.head = model.norm.clone(), quantised(model.head)

    def _run(self, tokens, mixer):
        stream = self.embed[tokens]
        h = torch.zeros(stream.shape, dtype=torch.bfloat16, device=stream.device)
        for i, m in enumerate(self.layers):
            q, scale, stream = cv.add_rmsnorm_int8(h, m["norm"], stream)
            w, ws, bias = m["proj_in"]
            x, forget, z = cv.int8_linear(q, scale, w, ws, bias).split(m["inner"], -1)
            q, scale = cv.quantize_int8(mixer(i, m, x, forget, z))
            w, ws, bias = m["proj_out"]
            h = cv.int8_linear(q, scale, w, ws, bias)
        q, scale, _ = cv.add_rmsnorm_int8(h, self.norm, stream)
        w, ws, _ = self.head
        return cv.int8_linear(q, scale, w, ws, out_dtype=torch.float32)

    @torch.no_grad()
    def prefill(self, tokens):
        """(logits, states): the prompt in one pass, one state per layer."""
        states = []

        def mixer(i, m, x, forget, z):
            y, state = cv.gated_linear_recurrence(x, forget, z, lower_bound=m["lower"])
            states.append(state)
            return y

        return self._run(tokens, mixer), states

    @torch.no_grad()
    def step(self, tokens, states):
        """Logits of one token per sequence; the states are updated in place."""
        return self._run(tokens, lambda i, m, x, forget, z: cv.gated_linear_recurrence_update(
            states[i], x, forget, z, lower_bound=m["lower"]))


def batch(batch_size, length, vocab, generator, motif=7):
    """Rows of two packed sequences, each a motif repeated; (tokens, reset)."""
    device = generator.device
    half = length // 2
    parts = []
    for n in (half, length - half):
        m = torch.randint(0, vocab, (batch_size, motif), device=device, generator=generator)
        parts.append(m.repeat(1, n // motif + 1)[:, :n])
    reset = torch.zeros(batch_size, length, dtype=torch.bool, device=device)
    reset[:, 0] = reset[:, half] = True
    return torch.cat(parts, 1), reset


def train(model, steps, generator, batch_size=32, length=129, vocab=64, lr=6e-3):
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        tokens, reset = batch(batch_size, length, vocab, generator)
        loss = F.cross_entropy(model(tokens[:, :-1], reset[:, :-1]).flatten(0, 1), tokens[:, 1:].flatten())
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return [float(v) for v in torch.stack(losses)]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--inner", type=int, default=768)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=64, help="tokens generated per sequence")
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    gen = torch.Generator(device="cuda").manual_seed(0)
    model = Model(width=args.width, inner=args.inner, layers=args.layers).cuda()
    losses = train(model, args.steps, gen)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} over {args.steps} steps")

    served = Served(model)
    prompt, _ = batch(8, 64, 64, gen)
    prompt = prompt[:, :32]
    with torch.no_grad():
        full = model(prompt)
    logits, states = served.prefill(prompt)
    off = float((logits - full).norm() / full.norm())
    print(f"int8 logits differ from the bfloat16 model's by {off:.3%} of their norm")

    token = logits[:, -1].argmax(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                 # a first step outside the graph, on copies of the states
        served.step(token, [s.clone() for s in states])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token.copy_(served.step(token, states).argmax(-1))
    out = [token.clone()]
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(args.tokens - 1):
        graph.replay()
        out.append(token.clone())
    torch.cuda.synchronize()
    each = (time.perf_counter() - began) / max(1, args.tokens - 1)
    check_errors()
    generated = torch.stack(out, 1)
    print(f"{each * 1e6:.0f} us a decode step of {len(prompt)} sequences, {args.layers} layers")
    return dict(losses=losses, off=off, prompt=prompt, generated=generated, served=served)


if __name__ == "__main__":
    main()
