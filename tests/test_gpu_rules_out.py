"""process_logits' out and autograd, on the GPU."""
import pytest
import torch

from sdmchat_amd import core

pytestmark = pytest.mark.gpu


def test_out_that_requires_a_gradient_is_refused():
    z = torch.randn(2, 50, device="cuda")
    out = torch.zeros(2, 50, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="inference"):
        core.process_logits(z, bias=torch.ones(50, device="cuda"), out=out)
    with torch.no_grad():
        core.process_logits(z, bias=torch.ones(50, device="cuda"), out=out)
    assert torch.equal(out.detach(), z + 1)


def test_a_graph_that_saved_the_logits_notices_that_they_were_overwritten():
    h = torch.randn(2, 50, device="cuda", requires_grad=True)
    z = h * 2
    loss = (z * z).sum()   # saves z
    core.process_logits(z.detach(), bias=torch.ones(50, device="cuda"), out=z.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors():
    with torch.inference_mode():
        z = torch.randn(2, 50, device="cuda")
        want = z + 1
        assert torch.equal(core.process_logits(z, bias=torch.ones(50, device="cuda"), out=z), want)


def test_logits_shared_by_another_allocation_record():
    """A tensor that shares the logits' memory without sharing their storage object (through dlpack) overlaps all the same."""
    z = torch.randn(6, 50, device="cuda")
    other = torch.utils.dlpack.from_dlpack(torch.utils.dlpack.to_dlpack(z[1:]))
    with pytest.raises(ValueError, match="overlaps"):
        core.process_logits(z[:5], bias=torch.ones(50, device="cuda"), out=other)
