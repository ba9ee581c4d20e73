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
