"""Host-side checks of the language-model operators' C structs (no GPU): the ctypes
mirrors equal what a C compiler makes of the header, field by field, and every op
has a status word."""

import ctypes
import pathlib
import re
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "ssm_b200.h"


def _structs():
    from metal_kernelops_b200 import _native as nat
    return (("ssm_add_rmsnorm_params", nat.AddRmsNormParams),
            ("ssm_int8_linear_params", nat.Int8LinearParams),
            ("ssm_gated_recurrence_params", nat.GatedRecurrenceParams),
            ("ssm_gated_recurrence_step_params", nat.GatedRecurrenceStepParams))


def test_fields_match_the_header():
    text = HEADER.read_text()
    for cname, struct in _structs():
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for decl in body.split(";"):
            decl = decl.strip()
            if decl:
                names = decl.split(None, 1)[1] if not decl.startswith("const") else decl.split(None, 2)[2]
                fields += [n.strip().lstrip("*").strip() for n in names.split(",")]
        assert [f for f, _ in struct._fields_] == fields, cname


def test_offsets_match_the_c_compiler(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include "ssm_b200.h"', "int main(void) {"]
    want = []
    for cname, struct in _structs():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(struct))
        for name, _ in struct._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {name}));')
            want.append(getattr(struct, name).offset)
    lines += ["return 0;", "}"]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines))
    subprocess.run([gcc, "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def test_status_words():
    from metal_kernelops_b200 import _native as nat
    assert {"add_rmsnorm", "int8_linear", "gated_recurrence"} <= set(nat.STATUS_SLOTS)
    assert nat.STATUS_SLOTS.index("selftest") == 7          # the words that were there keep their places


def test_oracle_definitions():
    """The 64-bit definitions against a second form of themselves: the recurrence's
    closed sum over the past, the norm's scale invariance, exact integer products."""
    import torch
    from oracle import lm_oracle as lm
    g = torch.Generator().manual_seed(0)
    x, f = (torch.randn(1, 9, 3, generator=g, dtype=torch.float64) for _ in range(2))
    low = torch.rand(3, generator=g, dtype=torch.float64)
    h0 = torch.randn(1, 3, generator=g, dtype=torch.float64)
    y, last = lm.gated_recurrence_ref(x, f, None, low, h0)
    keep = low + (1 - low) * torch.sigmoid(f)
    for t in range(9):
        want = h0 * keep[:, :t + 1].prod(1)
        for s in range(t + 1):
            want = want + keep[:, s + 1:t + 1].prod(1) * (1 - keep[:, s]) * x[:, s]
        torch.testing.assert_close(y[:, t], want, rtol=1e-12, atol=1e-12)
    assert torch.equal(last, y[:, -1])
    v, w = torch.randn(4, 16, generator=g, dtype=torch.float64), torch.ones(16, dtype=torch.float64)
    a, _ = lm.add_rmsnorm_ref(v, w, eps=0.0)
    b, _ = lm.add_rmsnorm_ref(v * 7, w, eps=0.0)
    torch.testing.assert_close(a, b, rtol=1e-13, atol=1e-13)
    q = torch.randint(-127, 128, (3, 20), generator=g, dtype=torch.int8)
    one = torch.ones(3)
    assert torch.equal(lm.int8_linear_ref(q, one, q, one).long(), q.long() @ q.long().t())


def test_norm_gradient_formula_against_autograd():
    import torch
    from oracle import lm_oracle as lm
    g = torch.Generator().manual_seed(1)
    x, res, dy, ds = (torch.randn(5, 12, generator=g, dtype=torch.float64) for _ in range(4))
    w = torch.randn(12, generator=g, dtype=torch.float64)
    for t in (x, res, w):
        t.requires_grad_(True)
    s = x + res
    y = w * s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    dx, dr, dw = torch.autograd.grad((y, s), (x, res, w), (dy, ds))
    d, dwf = lm.add_rmsnorm_grads_ref(dy, ds, s.detach(), w.detach())
    torch.testing.assert_close(d, dx)
    torch.testing.assert_close(d, dr)
    torch.testing.assert_close(dwf, dw)
