"""The distillation loss and its gradient through the C interface, loss and gradient in calls of their own, against float64
(tolerances: tests/test_gpu_distill.py)."""
import ctypes

import pytest
import torch

from sdmchat_amd import _lib, core
from tests._gpu_util import say
from tests.test_gpu_distill import U, make, reference

pytestmark = pytest.mark.gpu
REDUCTIONS = {"none": _lib.SDM_RT_NONE, "mean": _lib.SDM_RT_MEAN, "sum": _lib.SDM_RT_SUM}


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("N,V,K,dtype", [(1, 50, 3, torch.float32), (40, 1003, 12, torch.float32), (300, 2049, 5, torch.bfloat16),
                                         (5, 70001, 30, torch.bfloat16)])
def test_loss_then_gradient(reduction, along, N, V, K, dtype):
    """stats carry all that sdm_rt_distill_grad needs, whether or not the loss made a gradient along with itself."""
    say(f"[distill abi] {reduction} along={along} N={N} V={V} K={K} {dtype}")
    tau, alpha, lib = 1.5, 0.6, _lib.load()
    z, ids, top, lab = make(N, V, K, dtype, N + V)
    zd, idd, td, ld = z.cuda(), ids.cuda(), top.cuda(), lab.cuda()
    dims = _lib.SdmRtDistill(N, V, K, tau, alpha, -100, REDUCTIONS[reduction])
    head = (ctypes.byref(dims), zd.data_ptr(), V, core._DT[dtype], idd.data_ptr(), K, td.data_ptr(), K, ld.data_ptr())
    nbytes = lib.sdm_rt_distill_workspace_bytes(ctypes.byref(dims))
    ws = torch.empty(nbytes // 8 + 1, dtype=torch.long, device="cuda")
    loss = torch.empty(N if reduction == "none" else 1, device="cuda")
    stats = torch.full((N, 4), float("nan"), device="cuda")
    dz, first = torch.empty_like(zd), torch.empty_like(zd)
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.sdm_rt_distill_loss(*head, loss.data_ptr(), stats.data_ptr(), first.data_ptr() if along else None, V,
                                       ws.data_ptr(), nbytes, st))
    go = torch.full((N if reduction == "none" else 1,), 0.7, device="cuda")
    _lib.check(lib.sdm_rt_distill_grad(*head, stats.data_ptr(), go.data_ptr(), 0, dz.data_ptr(), V, st))
    rows, grad, lb, gb, target, n = reference(z, ids, top, lab, tau, alpha, reduction, grad_out=go.cpu())
    s = 1.0 / n if reduction == "mean" else 1.0
    if reduction == "none":
        assert bool(((loss.double().cpu() - rows).abs() <= lb).all())
    else:
        want = float(rows.sum()) * s
        assert abs(float(loss) - want) <= float(lb[target].sum()) * s + 2 * U * abs(want) + 1e-45
    half = torch.finfo(dtype).eps / 2
    err = (dz.double().cpu() - grad).abs()
    assert bool((err <= gb * (1 + half) + half * grad.abs() + 2.0 ** -126).all())
    assert not dz.cpu()[~target].any()
    if along:   # the gradient for an outer one of 1 (of the losses' sum for "none")
        err = (first.double().cpu() * 0.7 - grad).abs()
        # 0.7 times a rounded value, against the value for float32's 0.7 (off by 2^-25 of it)
        assert bool((err <= gb * (1 + half) + (half + U) * grad.abs() + 2.0 ** -126).all())


def _setup(seed=31):
    z, ids, top, lab = make(20, 700, 6, torch.float32, seed)
    return z, ids, top, lab, tuple(t.cuda() for t in (z, ids, top, lab))


def _want(z, ids, top, lab, go):
    _, grad, _, gb, _, _ = reference(z, ids, top, lab, 2.0, 0.5, grad_out=torch.tensor(go))
    return grad, gb + U * grad.abs() + 2.0 ** -126


def test_a_backward_captured_alone_replays_whatever_became_of_its_gradient():
    """The loss eager, its backward in a graph: every replay gives the gradient for what comes in then, also where the caller
    has written into the last one."""
    z, ids, top, lab, (zd, idd, td, ld) = _setup()
    go, stream = torch.ones((), device="cuda"), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        zz = zd.detach().requires_grad_(True)
        loss = core.distill_loss(zz, idd, td, labels=ld, alpha=0.5, temperature=2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        dz, = torch.autograd.grad(loss, zz, go, retain_graph=True)
    for x in (1.0, 3.0, 1.0, 0.0, 1.0):
        go.fill_(x)
        graph.replay()
        torch.cuda.synchronize()
        want, tol = _want(z, ids, top, lab, x)
        assert bool(((dz.double().cpu() - want).abs() <= tol).all()), x
        dz.fill_(5.0)   # the caller owns it between the replays
    with torch.cuda.stream(stream):   # the graph of the eager loss is whole
        eager, = torch.autograd.grad(loss, zz, torch.ones((), device="cuda"))
    torch.cuda.synchronize()
    want, tol = _want(z, ids, top, lab, 1.0)
    assert bool(((eager.double().cpu() - want).abs() <= tol).all())


def test_loss_and_backward_in_graphs_of_their_own():
    """Two backward replays after one of the loss, with other gradients coming in and the last result overwritten."""
    z, ids, top, lab, (zd, idd, td, ld) = _setup(32)
    go, stream = torch.ones((), device="cuda"), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    args = dict(labels=ld, alpha=0.5, temperature=2.0)
    with torch.cuda.stream(stream):
        zz = zd.detach().requires_grad_(True)
        torch.autograd.grad(core.distill_loss(zz, idd, td, **args), zz, go)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=stream):
        loss = core.distill_loss(zz, idd, td, **args)
    with torch.cuda.graph(second, stream=stream, pool=first.pool()):
        dz, = torch.autograd.grad(loss, zz, go, retain_graph=True)
    for r in range(3):
        z, ids, top, lab = make(20, 700, 6, torch.float32, 40 + r)
        for old, new in zip((zd, idd, td, ld), (z, ids, top, lab)):
            old.copy_(new)
        first.replay()
        for x in (1.0, -2.0, 1.0):
            go.fill_(x)
            second.replay()
            torch.cuda.synchronize()
            want, tol = _want(z, ids, top, lab, x)
            assert bool(((dz.double().cpu() - want).abs() <= tol).all()), (r, x)
            dz.zero_()
