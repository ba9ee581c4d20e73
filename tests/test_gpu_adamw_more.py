"""More of core.adamw and the AdamW optimiser on the GPU (test_gpu_adamw.py has the formula's twin and the bounds)."""
import io

import pytest
import torch

from sdmchat_amd import AdamW
from tests.test_gpu_adamw import SIZES, regrad, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_read_on_the_cpu_with_a_rate_on_the_device(bits):
    """The optimiser goes on where the saved one was, its schedule's tensor reaches it, also in a step captured after."""
    ps, gs = tensors(SIZES, [torch.float32, torch.bfloat16], 21)

    def fresh():
        qs = [torch.nn.Parameter(p.clone()) for p in ps]
        rate = torch.full((), 1e-3, device="cuda")
        return qs, rate, AdamW([dict(params=qs[:4]), dict(params=qs[4:])], lr=rate, state_bits=bits, capturable=True, seed=3)

    def give(qs, seed):
        for q, g in zip(qs, regrad(gs, seed)):
            if q.grad is None:
                q.grad = g
            else:
                q.grad.copy_(g)
    a, rate_a, oa = fresh()
    for s in range(3):
        give(a, s)
        rate_a.fill_(1e-3 * (s + 1))
        oa.step()
    f = io.BytesIO()
    torch.save(dict(p=[q.detach() for q in a], o=oa.state_dict()), f)
    f.seek(0)
    blob = torch.load(f, weights_only=True, map_location="cpu")
    b, rate_b, ob = fresh()
    with torch.no_grad():
        for q, v in zip(b, blob["p"]):
            q.copy_(v)
    ob.load_state_dict(blob["o"])
    assert torch.equal(rate_a, rate_b) and all(g["lr"] is rate_b for g in ob.param_groups)

    def same():
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(v, ob.state[y][k]) for x, y in zip(a, b) for k, v in oa.state[x].items())
    for s in range(3, 5):
        for qs, rate, opt in ((a, rate_a, oa), (b, rate_b, ob)):
            give(qs, s)
            rate.fill_(2e-3 * s)
            opt.step()
        same()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for s in range(5, 8):
        for qs, rate in ((a, rate_a), (b, rate_b)):
            give(qs, s)
            rate.fill_(1e-3 * s)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        same()
