"""int8_linear from several host threads at once: calls of one kernel with different numbers of
shared-memory stages do not refuse one another's launches, and their results stay right."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _call(tokens, k, features, seed):
    """A prepared call of the C entry, so that the threads spend their time in it, and its tensors."""
    from metal_kernelops_b200 import _native as nat
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-1, 2, (tokens, k), device="cuda", dtype=torch.int8, generator=g)
    w = torch.randint(-1, 2, (features, k), device="cuda", dtype=torch.int8, generator=g)
    xs, ws = torch.ones(tokens, device="cuda"), torch.ones(features, device="cuda")
    out = torch.empty(tokens, features, device="cuda")
    stream = torch.cuda.Stream()
    p = nat.Int8LinearParams(tokens, k, features, 0, 0, nat.SSM_F32, 0, x.data_ptr(), xs.data_ptr(), w.data_ptr(),
                             ws.data_ptr(), None, out.data_ptr(), None, 0, nat.status_word(x.device, "int8_linear"))
    return p, out, stream, (x, w, xs, ws)


@pytest.mark.parametrize("tokens", [1, 100])
def test_threads_with_different_shapes(tokens):
    from metal_kernelops_b200 import _native as nat
    lib = nat.lib()
    calls = [_call(tokens, k, 128, i) for i, k in enumerate((16384, 256, 16384, 512, 256, 8192))]
    torch.cuda.synchronize()
    refused, go = [], threading.Barrier(len(calls))

    def work(p, stream):
        torch.cuda.set_device(0)
        go.wait()
        for i in range(4000):
            if lib.ssm_int8_linear_fwd(p, stream.cuda_stream) != nat.SSM_OK:
                refused.append(lib.ssm_last_error())
            if i % 500 == 499:
                stream.synchronize()

    threads = [threading.Thread(target=work, args=(p, stream)) for p, _, stream, _ in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, (len(refused), refused[0])
    for _, out, _, (x, w, _, _) in calls:
        assert torch.equal(out, x.float() @ w.float().t())
