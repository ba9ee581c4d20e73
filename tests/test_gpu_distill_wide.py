"""The distillation loss's other kernels at sizes where their loops go round: the gradient from kept maxima and sums ("none",
and any gradient but 1 coming in), over several pieces of a thread and more rows than workgroups, and the loss without a
gradient, over several chunks of a row.  Against float64, tolerances as in tests/test_gpu_distill.py."""
import pytest
import torch

from sdmchat_amd import core
from tests._gpu_util import say
from tests.test_gpu_distill import U, check, make, reference

pytestmark = pytest.mark.gpu


def _repeat(ids, top):
    """Every other row names ids twice, one row one id throughout."""
    K = ids.shape[1]
    if K > 1:
        ids[::2, K // 2:] = ids[::2, :K - K // 2]
    ids[-1] = 11
    return ids, top


SHAPES = [(12, 4099, 9, 1.0, 0.4), (9, 4099, 1024, 1.5, 0.5), (10, 32003, 50, 2.0, 0.5), (7, 32003, 200, 1.0, 1.0),
          (6, 65541, 64, 1.5, 0.3), (5, 151936, 100, 2.0, 0.9), (5, 151936, 20, 1.5, 0.5), (4, 300001, 33, 1.0, 0.5),
          (3, 300001, 7, 2.5, 0.6)]


@pytest.mark.parametrize("N,V,K,tau,alpha", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_gradient_from_kept_sums(N, V, K, tau, alpha, dtype, reduction):
    say(f"[distill grad] {reduction} N={N} V={V} K={K} tau={tau} alpha={alpha} {dtype}")
    z, ids, top, lab = make(N, V, K, dtype, N + V + K + 1, labels=alpha < 1, empty=False)
    ids, top = _repeat(ids, top)
    if lab is not None:
        lab[::3] = ids[::3, 0]
        lab[1] = -100
    ids[2] = -1
    go = torch.linspace(-1.5, 2.0, N) if reduction == "none" else torch.tensor(0.3)
    check(z, ids, top, lab, tau, alpha, reduction, grad_out=go)


@pytest.mark.parametrize("N,V,K,tau,dtype", [(2700, 1003, 9, 2.0, torch.float32), (1300, 4099, 5, 1.5, torch.bfloat16),
                                             (1025, 2049, 70, 1.0, torch.float32), (66000, 37, 3, 1.5, torch.float32)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_more_rows_than_workgroups(N, V, K, tau, dtype, reduction):
    """A workgroup takes several rows in turn, with and without a target, repeated ids among them."""
    z, ids, top, lab = make(N, V, K, dtype, N, empty=False)
    ids, top = _repeat(ids, top)
    gone = torch.rand(N, generator=torch.Generator().manual_seed(3)) < 0.2
    ids[gone], lab[gone] = -1, -100
    z[gone] = float("nan")
    go = torch.linspace(-1.5, 2.0, N) if reduction == "none" else torch.tensor(0.3)
    check(z, ids, top, lab, tau, 0.5, reduction, grad_out=go)


@pytest.mark.parametrize("N,V,K,tau,alpha", SHAPES + [(700, 2049, 9, 1.0, 0.5), (3, 600001, 5, 1.0, 0.5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_alone(N, V, K, tau, alpha, dtype):
    """No gradient recorded: rows in chunks, their largest value in the first, a middle or the last one or in the tail, rows
    that rise all along, and rows that begin with -inf."""
    z, ids, top, lab = make(N, V, K, dtype, N + V + K + 2, labels=alpha < 1)
    for r, at in ((0, 0), (1, V - 1), (2, V // 2)):
        z[r, at] = 40.0
    if N > 4:
        z[3] = torch.linspace(-60, 60, V).to(dtype)
        z[4, :V // 2] = float("-inf")
        ids[4] = torch.where(ids[4] >= 0, ids[4].clamp(min=V // 2), ids[4])   # a target that is not masked
        if lab is not None:
            lab[4] = V - 1
    args = dict(temperature=tau, labels=None if lab is None else lab.cuda(), alpha=alpha)
    rows, _, lb, _, target, n = reference(z, ids, top, lab, tau, alpha)
    with torch.no_grad():
        got = {r: core.distill_loss(z.cuda(), ids.cuda(), top.cuda(), reduction=r, **args).double().cpu() for r in ("none", "mean", "sum")}
    assert bool(((got["none"] - rows).abs() <= lb).all())
    want, tol = float(rows.sum()), float(lb[target].sum())
    assert abs(float(got["sum"]) - want) <= tol + 2 * U * abs(want)
    assert abs(float(got["mean"]) - want / n) <= tol / n + 2 * U * abs(want) / n
