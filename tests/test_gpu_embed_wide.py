"""The embedding's gradient on both sides of the width that one launch takes, against float64 (tolerances:
tests/test_gpu_embed.py)."""
import pytest
import torch

from sdmchat_amd import core
from tests.test_gpu_embed import _check_grad, _ids

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [1021, 1024, 1025, 1032, 2050, 4096])
@pytest.mark.parametrize("N", [1, 63, 700, 5120])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widths_around_one_launch(d, N, dtype):
    g = torch.Generator().manual_seed(N + d)
    for kind in ("zipf", "one", "bytes"):
        ids = _ids(kind, N, 600, g)
        pad = None if kind == "one" else int(ids[-1])
        dy = torch.randn(N, d, generator=g).to(dtype)
        got = core.embedding_backward(ids.cuda(), dy.cuda(), 600, 1.3, pad)
        _check_grad(got, ids, dy, 600, 1.3, pad)
        assert torch.equal(got, core.embedding_backward(ids.cuda(), dy.cuda(), 600, 1.3, pad))
