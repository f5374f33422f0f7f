"""The operators together: the example model trains, and its int8 form serves.

Checked: training lowers the loss below what guessing gives; a gradient step equals
the 64-bit model's (the operators' definitions in ``oracle.lm_oracle``); the int8
logits stay near the trained model's; prefill and token-by-token decoding agree; the
captured decode step generates what stepping by hand does.
"""

import importlib.util
import math
import pathlib

import pytest
import torch
import torch.nn.functional as F

from oracle import lm_oracle as lm

pytestmark = pytest.mark.gpu


def _example():
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "recurrent_lm.py"
    spec = importlib.util.spec_from_file_location("recurrent_lm", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_trains_and_serves():
    ex = _example()
    got = ex.main(["--layers", "2", "--width", "128", "--inner", "200", "--steps", "80", "--tokens", "12"])
    assert got["losses"][-1] < 0.7 * math.log(64) < got["losses"][0]
    # two quantisations of half a step in 127 per product, over two layers and the head
    assert got["off"] < 0.1
    served, prompt, generated = got["served"], got["prompt"], got["generated"]
    # the captured steps against steps by hand from the same prompt
    logits, states = served.prefill(prompt)
    token = logits[:, -1].argmax(-1)
    for i in range(generated.shape[1]):
        assert torch.equal(token, generated[:, i])
        token = served.step(token, states).argmax(-1)
    # decoding the prompt token by token from empty states against one pass over it
    whole, final = served.prefill(prompt)
    states = [torch.zeros_like(s) for s in final]
    steps = torch.stack([served.step(prompt[:, i], states) for i in range(prompt.shape[1])], 1)
    # the same operations on rows alike; a state's last bits may move a bf16 rounding or a quantised value by a step
    assert float((steps - whole).norm() / whole.norm()) < 2e-2
    for a, b in zip(states, final):
        assert float((a - b).norm() / b.norm()) < 2e-2


def test_gradients_equal_the_definition():
    """One packed batch through the bf16 model against float64, norm-relative 3e-2:
    bf16 activations (2^-8 each) through a handful of products."""
    ex = _example()
    torch.manual_seed(1)
    model = ex.Model(vocab=16, width=64, inner=48, layers=2).cuda()
    gen = torch.Generator(device="cuda").manual_seed(2)
    tokens, reset = ex.batch(3, 41, 16, gen)
    loss = F.cross_entropy(model(tokens[:, :-1], reset[:, :-1]).flatten(0, 1), tokens[:, 1:].flatten())
    loss.backward()
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in model.named_parameters()}
    t, r = tokens.cpu(), reset.cpu()[:, :-1]
    stream = p["embed.weight"][t[:, :-1]]
    h = torch.zeros_like(stream)

    def norm(s, w):
        return w * s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)

    for i in range(2):
        stream = stream + h
        y = norm(stream, p[f"layers.{i}.norm"])
        proj = F.linear(y, p[f"layers.{i}.in_proj.weight"], p[f"layers.{i}.in_proj.bias"])
        x, forget, z = proj.split(48, -1)
        y, _ = lm.gated_recurrence_ref(x, forget, z, p[f"layers.{i}.lower"].clamp(0, 0.99), None, r)
        h = F.linear(y, p[f"layers.{i}.out_proj.weight"], p[f"layers.{i}.out_proj.bias"])
    logits = F.linear(norm(stream + h, p["norm"]), p["head.weight"])
    ref = F.cross_entropy(logits.flatten(0, 1), t[:, 1:].flatten())
    ref.backward()
    assert abs(float(loss.detach()) - float(ref.detach())) <= 2e-2 * float(ref.detach())
    for k, v in model.named_parameters():
        err = float((v.grad.double().cpu() - p[k].grad).norm() / (p[k].grad.norm() + 1e-12))
        assert err <= 3e-2, (k, err)
