"""The embedding under autograd's other modes, on the GPU."""
import pytest
import torch

from sdmchat_amd import core

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("needs", [False, True])
def test_a_tangent_is_refused(needs):
    """Forward-mode differentiation is not built: the tangent of a table is refused, not dropped."""
    ids, table = torch.tensor([1, 2, 2], device="cuda"), torch.randn(5, 8, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(table.clone().requires_grad_(needs), torch.ones_like(table))
        with pytest.raises(RuntimeError):
            core.embedding(ids, dual)
        assert torch.equal(core.embedding(ids, table, 2.0), table[ids] * 2.0)   # a table without one
    assert torch.equal(core.embedding(ids, table, 2.0), table[ids] * 2.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [700, 9000])
def test_a_recorded_gradient_is_the_kernels(dtype, N):
    """create_graph changes no bit of the gradient, which is the same from call to call."""
    g = torch.Generator().manual_seed(N)
    ids = torch.randint(0, 40, (N,), generator=g).cuda()
    table = torch.randn(300, 70, generator=g).to(dtype).cuda().requires_grad_(True)
    dy = torch.randn(N, 70, generator=g).to(dtype).cuda()

    def grad(again):
        return torch.autograd.grad(core.embedding(ids, table, 1.7, 3), table, dy, create_graph=again)[0].detach()
    want = grad(False)
    for _ in range(3):
        assert torch.equal(grad(True), want)


@pytest.mark.parametrize("pad", [None, 4])
def test_differentiated_twice_and_three_times(pad):
    """Gradients of gradients through the lookup, against torch's own embedding in float64: sums of 60 products each, three
    deep, each off by 2^-24 of its largest."""
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 9, (5, 12), generator=g).cuda()
    table, w = torch.randn(9, 6, generator=g).cuda(), torch.randn(5, 12, 6, generator=g).cuda()

    def chain(t, w, f):
        gr, = torch.autograd.grad((f(t) ** 3 * w).sum(), t, create_graph=True)
        g2, = torch.autograd.grad((gr ** 2).sum(), t, create_graph=True)
        g3, = torch.autograd.grad((g2 * t).sum(), t)
        return gr.detach(), g2.detach(), g3
    got = chain(table.clone().requires_grad_(True), w, lambda t: core.embedding(ids, t, 1.5, pad))
    want = chain(table.double().requires_grad_(True), w.double(), lambda t: torch.nn.functional.embedding(ids, t, pad) * 1.5)
    for a, b in zip(got, want):
        assert float((a - b).abs().max()) <= 3 * 64 * 2.0 ** -24 * float(b.abs().max()) * 4


def test_an_outer_gradient_that_is_expanded():
    """The rows that come into the second derivative may be one row repeated, or not contiguous."""
    ids = torch.tensor([0, 2, 2, 3], device="cuda")
    table = torch.randn(4, 6, device="cuda", requires_grad=True)
    dy = torch.randn(4, 6, device="cuda", requires_grad=True)
    gr, = torch.autograd.grad(core.embedding(ids, table, 2.0), table, dy, create_graph=True)
    for outer in (torch.ones(1, 1, device="cuda").expand(4, 6), torch.randn(6, 4, device="cuda").t()):
        got, = torch.autograd.grad(gr, dy, outer, retain_graph=True)
        assert torch.equal(got, outer[ids] * 2.0)
