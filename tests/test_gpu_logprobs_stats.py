"""sdm_rt_token_logprobs_grad on the statistics of a call that asked for no entropy: the log probabilities' gradient is theirs, the
entropy's is NaN rather than wrong."""
import ctypes

import pytest
import torch

from sdmchat_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [50, 5000, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 4])
def test_statistics_without_entropy(V, dtype, k):
    lib, N = _lib.load(), 5
    gen = torch.Generator().manual_seed(V + k)
    z = torch.randn(N, V, generator=gen).to(dtype).cuda()
    z[3] = -torch.inf
    y = torch.randint(0, V, (N,), generator=gen).cuda()
    y[4] = -100
    code = 0 if dtype == torch.float32 else 1
    dims = _lib.SdmRtLogprob(N, V, k, 0.9, -100)
    at = ctypes.byref(dims)
    nbytes = lib.sdm_rt_token_logprobs_workspace_bytes(at, code)
    ws = torch.empty(max(nbytes, 8), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    ids, tops = torch.empty(N, max(k, 1), dtype=torch.int64, device="cuda"), torch.empty(N, max(k, 1), device="cuda")
    g = torch.randn(N, generator=gen).cuda()

    def stats(entropy):
        lp, h, s = torch.empty(N, device="cuda"), torch.empty(N, device="cuda"), torch.empty(N, 4, device="cuda")
        _lib.check(lib.sdm_rt_token_logprobs(at, z.data_ptr(), V, code, y.data_ptr(), lp.data_ptr(), h.data_ptr() if entropy else None,
                                             ids.data_ptr(), tops.data_ptr(), s.data_ptr(), ws.data_ptr(), nbytes, stream))
        return s

    def grad(s, dlp, dh):
        dz = torch.empty_like(z)
        _lib.check(lib.sdm_rt_token_logprobs_grad(at, z.data_ptr(), V, code, y.data_ptr(), s.data_ptr(), dlp, 1, dh, 1, dz.data_ptr(), V,
                                                  stream))
        return dz
    with_h, without = stats(True), stats(False)
    assert torch.equal(with_h[:, :2], without[:, :2])
    want = grad(with_h, g.data_ptr(), None)
    assert torch.equal(grad(without, g.data_ptr(), None), want) and bool(want[0].any()) and not want.isnan().any()
    assert not want[3:].any()   # a row of -inf, a row without a target
    assert not grad(with_h, g.data_ptr(), g.data_ptr()).isnan().any()
    for dlp in (None, g.data_ptr()):
        bad = grad(without, dlp, g.data_ptr())
        assert bool(bad[[0, 1, 2, 4]].isnan().all()) and not bad[3].any()
    zero = torch.zeros_like(g)
    assert not grad(without, None, zero.data_ptr()).any()
