"""core.token_logprobs where a slice lists more keys than are ranked at once (over 2 top + 64): one wave narrows the list while
the others go on to the next barrier.  Many rows of many waves in one call, against the definitions."""
import pytest
import torch

from sdmchat_amd import core
from tests.test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


def rows(N, V, dtype, k, seed):
    """Logits whose greatest lie in the 16-byte pieces of a few threads, several of them a thread, all different where the type
    allows; each row has its own threads and its own number of them."""
    g = torch.Generator().manual_seed(seed)
    kn = 8 if dtype == torch.bfloat16 else 4
    z = torch.randn(N, V, generator=g)
    for r in range(N):
        pieces = torch.randperm(V // kn, generator=g)[:k + 1 + r % (k // 2 + 8)]
        at = (pieces[:, None] * kn + torch.arange(kn)).reshape(-1)
        z[r, at] = 8.0 + 4.0 * torch.rand(len(at), generator=g)
    return z.to(dtype), torch.randint(0, V, (N,), generator=g)


@pytest.mark.parametrize("V", [4096, 32768, 32003, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [3, 30, 100])
def test_lists_that_are_narrowed(V, dtype, k):
    z, y = rows(48, V, dtype, k, V + k)
    check(z, y, 1.0, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_lists_in_many_workgroups_at_once(dtype):
    """Workgroups of every kind side by side, several to a compute unit: each row's alternatives are those of its first copy."""
    k, copies = 64, 40
    z, _ = rows(32, 32768, dtype, k, 7)
    z[::4] = torch.randn(8, 32768, generator=torch.Generator().manual_seed(8)).to(dtype)   # rows without a long list
    z[1::8] = (z[1::8].float() * 0.5).round().to(dtype)   # and rows of ties
    one = core.token_logprobs(z.cuda(), None, top=k)
    want = torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(one.top_ids.cpu(), want)
    many = core.token_logprobs(z.cuda().repeat(copies, 1), None, top=k)
    assert torch.equal(many.top_ids, one.top_ids.repeat(copies, 1))
    assert torch.equal(many.top_logprobs, one.top_logprobs.repeat(copies, 1))
