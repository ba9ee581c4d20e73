"""core.distill_loss and its gradient on the GPU against the definitions in float64.

Tolerances, per row, with A the largest |z - max| / min(temperature, 1) and c the length of a thread's chain of sums: an
exponential is off by at most (1 + A) 2^-23 relative (two float32 roundings of its argument and the unit's own last place),
a sum of them by c 2^-24 more, so p by rel = 2^-24 (c + 4 (2 + A)).  A row's loss is a weighted mean of log-probabilities
of size up to A + log(vocab), off by rel + 2^-22 (A + 12); a gradient by rel of each of its terms and the last rounding
(eps / 2)."""
import math

import pytest
import torch

from sdmchat_amd import OneSdmLM, core
from tests._gpu_util import say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(N, V, K, dtype, seed, labels=True, spread=3.0, empty=True):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(N, V, generator=g) * spread).to(dtype)
    ids = torch.randint(0, V, (N, K), generator=g)
    top = torch.randn(N, K, generator=g) * 2
    lab = torch.randint(0, V, (N,), generator=g) if labels else None
    if empty and N > 4:
        ids[1] = -1
        if K:
            ids[2, K // 2:] = -1
            ids[3, 0] = V + 5
        if labels:
            lab[0] = -100
            lab[1] = -100
    return z, ids, top, lab


def reference(z, ids, top, lab, tau, alpha, reduction="mean", ignore=-100, grad_out=None):
    """Losses, gradient, and the per-row bounds of their errors, in float64 on the CPU."""
    N, V = z.shape
    z = z.double()
    live = (ids >= 0) & (ids < V) & (top.double() / tau > -math.inf) & (alpha > 0)
    has_t = live.any(1) if ids.shape[1] else torch.zeros(N, dtype=torch.bool)
    t = torch.where(live, top.double() / tau, -math.inf)
    q = torch.softmax(t, 1) if ids.shape[1] else t
    q = torch.where(live, q, 0.0)
    logp = torch.log_softmax(z / tau, 1)
    at = ids.clamp(0, V - 1)
    terms = torch.where(q > 0, q * (torch.log(q) - logp.gather(1, at)), torch.where(q != q, q, 0.0))
    loss = torch.where(has_t, alpha * tau ** 2 * terms.sum(1), 0.0)
    grad = torch.where(has_t[:, None], alpha * tau * (logp.exp() - torch.zeros_like(z).scatter_add(1, at, q)), 0.0)
    size = torch.where(has_t[:, None], alpha * tau * (logp.exp() + torch.zeros_like(z).scatter_add(1, at, q)), 0.0)
    has_y = torch.zeros(N, dtype=torch.bool)
    if lab is not None and alpha < 1:
        has_y = (lab >= 0) & (lab < V) & (lab != ignore)
        y = lab.clamp(0, V - 1)[:, None]
        lp1 = torch.log_softmax(z, 1)
        loss = loss + torch.where(has_y, -(1 - alpha) * lp1.gather(1, y)[:, 0], 0.0)
        hot = torch.zeros_like(z).scatter(1, y, 1.0)
        grad = grad + torch.where(has_y[:, None], (1 - alpha) * (lp1.exp() - hot), 0.0)
        size = size + torch.where(has_y[:, None], (1 - alpha) * (lp1.exp() + hot), 0.0)
    target = has_t | has_y
    n = max(int(target.sum()), 1)
    w = torch.full((N,), 1.0 / n if reduction == "mean" else 1.0, dtype=torch.float64) * target
    if grad_out is not None:
        w = w * grad_out.double()
    finite = torch.where(z.isfinite(), z, 0.0)
    A = ((finite.amax(1) - finite.amin(1)) / min(tau, 1.0)).clamp(max=150.0)   # below exp(-150) a term is nothing
    rel = U * (V / 64 + 16 + 4 * (2 + A))
    lbound = (alpha * tau ** 2 + 1) * (rel + 4 * U * (A + 12)) + 4 * U * loss.abs()
    gbound = rel[:, None] * size * w.abs()[:, None]
    return loss, grad * w[:, None], lbound, gbound, target, n


def check(z, ids, top, lab, tau, alpha, reduction="mean", ignore=-100, grad_out=None):
    z_d = z.cuda().requires_grad_(True)
    loss = core.distill_loss(z_d, ids.cuda(), top.cuda(), temperature=tau, labels=None if lab is None else lab.cuda(),
                             alpha=alpha, ignore_index=ignore, reduction=reduction)
    go = torch.ones_like(loss) if grad_out is None else grad_out.float().cuda().reshape(loss.shape)
    dz, = torch.autograd.grad(loss, z_d, go)
    rows, grad, lb, gb, target, n = reference(z, ids, top, lab, tau, alpha, reduction, ignore, grad_out)
    got = loss.detach().double().cpu()
    if reduction == "none":
        assert bool(((got - rows).abs() <= lb).all())
    else:
        s = 1.0 / n if reduction == "mean" else 1.0
        want = float(rows.sum()) * s
        assert abs(float(got) - want) <= float(lb[target].sum()) * s + 2 * U * abs(want) + 1e-45
    half = torch.finfo(z.dtype).eps / 2
    err = (dz.double().cpu() - grad).abs()
    # float32's smallest normal number is where the exponential unit ends
    tol = gb * (1 + half) + half * grad.abs() + 2.0 ** -126
    assert bool((err <= tol).all()), float((err - tol).max())
    assert not dz.cpu()[~target].any()
    return loss, dz


@pytest.mark.parametrize("N,V,K,tau,alpha", [
    (1, 1, 1, 1.0, 1.0), (1, 2, 1, 2.0, 0.5), (7, 5, 9, 1.0, 0.3), (6, 63, 3, 1.5, 1.0), (5, 64, 64, 1.0, 0.7),
    (9, 257, 16, 4.0, 0.5), (33, 1000, 50, 2.0, 0.9), (64, 2048, 1, 1.0, 0.5), (12, 4099, 1024, 2.0, 0.5), (8, 8193, 0, 1.0, 0.0),
    (300, 32768, 32, 2.0, 0.5), (40, 32003, 100, 1.0, 1.0), (6, 65541, 20, 1.0, 0.5), (5, 131072, 20, 3.0, 0.4),
    (6, 151936, 64, 1.0, 0.5), (3, 262147, 5, 2.0, 0.5), (2, 600001, 5, 1.0, 0.5),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_and_gradient(N, V, K, tau, alpha, dtype):
    say(f"[distill] N={N} V={V} K={K} tau={tau} alpha={alpha} {dtype}")
    check(*make(N, V, K, dtype, N + V + K, labels=alpha < 1), tau, alpha)


@pytest.mark.parametrize("N,V,K,dtype", [(530, 66001, 5, torch.bfloat16), (300, 100008, 70, torch.bfloat16),
                                         (300, 34005, 20, torch.float32)])
def test_rows_in_turn(N, V, K, dtype):
    """More rows than compute units, each too long for several workgroups to a unit: a workgroup takes rows in turn, some of
    them without a target and full of NaN."""
    z, ids, top, lab = make(N, V, K, dtype, N)
    gone = torch.rand(N, generator=torch.Generator().manual_seed(2)) < 0.2
    gone[-3:] = True
    ids[gone], lab[gone] = -1, -100
    z[gone] = float("nan")
    check(z, ids, top, lab, 2.0, 0.5)


@pytest.mark.parametrize("V,dtype", [(98305, torch.float32), (200003, torch.bfloat16), (300001, torch.float32)])
def test_many_targets_of_rows_in_chunks(V, dtype):
    """Rows that pass in chunks, the first of them partial, with entries in all of them and around their edges."""
    z, ids, top, lab = make(40, V, 1024, dtype, V, empty=False)
    kn = 16 // z.element_size()
    whole, chunk = V // kn * kn, 16 * 768 * kn
    edges = torch.tensor([e + o for e in range(whole % chunk, V, chunk) for o in range(-kn, kn)] + [0, whole - 1, V - 1])
    edges = edges[(edges >= 0) & (edges < V)].unique()
    ids[:, :len(edges)] = edges
    lab[:len(edges)] = edges[:len(lab)]
    check(z, ids, top, lab, 2.0, 0.5)


@pytest.mark.parametrize("K", [2, 63, 64, 65, 200, 1024])
def test_repeated_ids(K):
    """Ids that repeat, among few and many entries, with the label among them or not."""
    z, ids, top, lab = make(24, 3001, K, torch.float32, K, empty=False)
    ids[8:16, K // 2:] = ids[8:16, :K - K // 2]
    ids[16:20] = 7
    lab[::2] = ids[::2, 0]
    check(z, ids, top, lab, 1.5, 0.5)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("go", [1.0, 0.125, -3.3, 0.0])
def test_reductions_and_outer_gradients(reduction, go):
    z, ids, top, lab = make(40, 1003, 12, torch.float32, 5)
    g = torch.randn(40, generator=torch.Generator().manual_seed(1)).double() if reduction == "none" else torch.tensor(go).double()
    check(z, ids, top, lab, 2.0, 0.6, reduction, grad_out=g.float())


def test_leading_dimensions_and_types_of_the_targets():
    z, ids, top, lab = make(24, 500, 6, torch.bfloat16, 6)
    a = core.distill_loss(z.cuda(), ids.cuda(), top.cuda(), labels=lab.cuda(), alpha=0.5, reduction="none")
    b = core.distill_loss(z.view(2, 3, 4, 500).cuda(), ids.view(2, 3, 4, 6).int().cuda(), top.view(2, 3, 4, 6).cuda(),
                          labels=lab.view(2, 3, 4).int().cuda(), alpha=0.5, reduction="none")
    assert tuple(b.shape) == (2, 3, 4) and torch.equal(a, b.reshape(-1))
    one = core.distill_loss(z[0].cuda(), ids[0].cuda(), top[0].bfloat16().cuda())
    assert one.dim() == 0 and math.isfinite(float(one))


def test_a_row_without_a_target_counts_nothing_whatever_it_holds():
    z, ids, top, lab = make(8, 300, 4, torch.float32, 7)
    ids[5], lab[5] = -1, -100
    z[5] = float("nan")
    z[1, 3] = float("inf")
    loss, dz = check(z, ids, top, lab, 2.0, 0.5)
    assert math.isfinite(float(loss.detach()))


def test_nothing_has_a_target():
    z, ids, top, lab = make(8, 300, 4, torch.float32, 8)
    for reduction in ("mean", "sum", "none"):
        loss, dz = check(z, torch.full_like(ids, -1), top, torch.full_like(lab, -100), 1.0, 0.5, reduction)
        assert not loss.any() and not dz.any()
    z0 = torch.zeros(0, 300, device="cuda", requires_grad=True)
    loss = core.distill_loss(z0, ids[:0].cuda(), top[:0].cuda(), labels=lab[:0].cuda(), alpha=0.5)
    loss.backward()
    assert float(loss.detach()) == 0.0 and tuple(z0.grad.shape) == (0, 300)
    assert tuple(core.distill_loss(z0, ids[:0].cuda(), top[:0].cuda(), reduction="none").shape) == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_vocabulary_and_teacher_entries(dtype):
    """-inf and the type's lowest value among the logits, -inf among the teacher's, repeated ids."""
    z, ids, top, lab = make(16, 400, 8, dtype, 9)
    z[:, ::3] = float("-inf")
    z[:, 1::3] = torch.finfo(dtype).min
    ids = ids // 3 * 3 + 2   # the teacher's tokens are not masked
    ids = ids.clamp(max=398)
    lab = lab // 3 * 3 + 2
    lab[lab > 398] = 2
    top[:, 1::2] = float("-inf")
    top[4] = float("-inf")   # no teacher at all
    ids[6] = 5               # one id, eight times
    lab[6] = 5
    check(z, ids, top, lab, 1.5, 0.5)


def test_a_teacher_token_that_the_student_masks():
    z, ids, top, _ = make(8, 100, 4, torch.float32, 10, labels=False)
    z[0, ids[0, 0]] = float("-inf")
    z_d = z.cuda().requires_grad_(True)
    rows = core.distill_loss(z_d, ids.cuda(), top.cuda(), reduction="none")
    assert float(rows[0]) == float("inf") and bool(rows[1:].isfinite().all())
    dz, = torch.autograd.grad(rows.sum(), z_d)
    _, grad, _, gb, _, _ = reference(z, ids, top, None, 1.0, 1.0, "sum")
    assert bool(((dz.double().cpu() - grad).abs() <= gb + U * grad.abs() + 2.0 ** -126).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_and_infinity_reach_their_row_alone(bad):
    z, ids, top, lab = make(8, 100, 4, torch.float32, 11)
    z[5, 50] = bad
    top[6, 0] = bad
    z_d = z.cuda().requires_grad_(True)
    rows = core.distill_loss(z_d, ids.cuda(), top.cuda(), labels=lab.cuda(), alpha=0.5, reduction="none")
    dz, = torch.autograd.grad(rows.sum(), z_d)
    assert bool(rows[5].isnan()) and bool(rows[6].isnan())
    rest = [0, 1, 2, 3, 4, 7]
    assert bool(rows[rest].isfinite().all()) and bool(dz[rest].isfinite().all())
    assert bool(dz[5].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    z, ids, top, lab = make(10, 999, 6, dtype, 12)
    want = core.distill_loss(z.cuda(), ids.cuda(), top.cuda(), labels=lab.cuda(), alpha=0.5, temperature=2.0, reduction="none")
    wide = torch.randn(10, 1300).to(dtype).cuda()
    wide[:, 5:1004] = z.cuda()
    views = [wide[:, 5:1004], z.t().contiguous().cuda().t()]
    for v in views:
        got = core.distill_loss(v, ids.t().contiguous().cuda().t(), top.repeat(1, 2).cuda()[:, :6], labels=lab.cuda(), alpha=0.5,
                                temperature=2.0, reduction="none")
        assert torch.equal(got, want)
    leaf = wide.clone().requires_grad_(True)
    core.distill_loss(leaf[:, 5:1004], ids.cuda(), top.cuda(), labels=lab.cuda(), alpha=0.5, temperature=2.0).backward()
    z_d = z.cuda().requires_grad_(True)
    core.distill_loss(z_d, ids.cuda(), top.cuda(), labels=lab.cuda(), alpha=0.5, temperature=2.0).backward()
    assert torch.equal(leaf.grad[:, 5:1004], z_d.grad) and not leaf.grad[:, :5].any() and not leaf.grad[:, 1004:].any()
    row = z[:1].cuda().expand(10, 999)   # one row of logits for ten targets
    got = core.distill_loss(row, ids.cuda(), top.cuda(), reduction="none")
    assert torch.equal(got, core.distill_loss(row.contiguous(), ids.cuda(), top.cuda(), reduction="none"))


def test_gradient_against_differences():
    """The loss along random sign vectors u: the difference quotient at h is off by h^2 / 6 of the third derivative, at most
    alpha / tau + (1 - alpha) times 1 (the third cumulant of values of +-1), and by the losses' errors over h."""
    z, ids, top, lab = make(6, 40, 5, torch.float32, 13, spread=1.0)
    tau, alpha, h = 2.0, 0.5, 0.03
    z_d = z.cuda().requires_grad_(True)
    args = dict(temperature=tau, labels=lab.cuda(), alpha=alpha, reduction="sum")
    loss = core.distill_loss(z_d, ids.cuda(), top.cuda(), **args)
    dz, = torch.autograd.grad(loss, z_d)
    lb = float(reference(z, ids, top, lab, tau, alpha, "sum")[2].sum())
    for s in range(4):
        u = (torch.randint(0, 2, z.shape, generator=torch.Generator().manual_seed(s)) * 2 - 1).float()
        with torch.no_grad():
            up, down = (float(core.distill_loss((z + k * h * u).cuda(), ids.cuda(), top.cuda(), **args)) for k in (1, -1))
        got = float((dz.cpu().double() * u.double()).sum())
        # z + h u is rounded too: 2^-24 of 4 in each of 40 places of a row
        tol = h * h / 6 * 6 * (alpha / tau + 1 - alpha) + (lb + 6 * 8 * U) / h
        assert abs(got - (up - down) / (2 * h)) <= tol


def test_backward_twice_and_not_differentiable_again():
    z, ids, top, lab = make(20, 333, 5, torch.bfloat16, 14)
    z_d = z.cuda().requires_grad_(True)
    loss = core.distill_loss(z_d, ids.cuda(), top.cuda())
    a, = torch.autograd.grad(loss, z_d, retain_graph=True)
    keep = a.clone()
    a.fill_(7.0)   # the caller owns its gradient
    b, = torch.autograd.grad(loss, z_d, retain_graph=True)
    c, = torch.autograd.grad(loss, z_d, torch.tensor(4.0, device="cuda"))
    assert torch.equal(keep, b) and torch.equal(c, b * 4)
    g, = torch.autograd.grad(core.distill_loss(z_d, ids.cuda(), top.cuda()), z_d, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_no_gradient_asked_for():
    z, ids, top, lab = make(20, 333, 5, torch.float32, 15)
    with torch.no_grad():
        a = core.distill_loss(z.cuda().requires_grad_(True), ids.cuda(), top.cuda())
    assert not a.requires_grad
    b = core.distill_loss(z.cuda().requires_grad_(True), ids.cuda(), top.cuda().requires_grad_(True))
    assert torch.equal(a, b.detach())
    b.backward()


def test_no_gradient_is_computed_where_none_is_recorded():
    """Under no_grad logits that require a gradient cost no more memory than ones that do not."""
    z, ids, top, lab = (t.cuda() for t in make(64, 32768, 5, torch.bfloat16, 18))
    z.requires_grad_(True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        core.distill_loss(z, ids, top, labels=lab, alpha=0.5)
    assert torch.cuda.max_memory_allocated() - before < z.numel() * z.element_size()


def test_refusals():
    z, ids, top, lab = (t.cuda() for t in make(6, 50, 4, torch.float32, 16))
    for args, kw, text in (((z.half(), ids, top), {}, "float32 or bfloat16"), ((z, ids[:5], top[:5]), {}, "top_ids"),
                           ((z, ids, top[:, :3]), {}, "top_ids"), ((z, ids.float(), top), {}, "int64"),
                           ((z, ids, top.long()), {}, "floating"), ((z, ids, top), dict(labels=lab[:5], alpha=0.5), "labels"),
                           ((z, ids, top), dict(labels=lab.float(), alpha=0.5), "int64"), ((z, ids, top), dict(alpha=0.5), "alpha"),
                           ((z, ids, top), dict(reduction="max"), "reduction"), ((z, ids.cpu(), top), {}, "cpu"),
                           ((z[:, :0], ids, top), {}, "vocab")):
        with pytest.raises(ValueError, match=text):
            core.distill_loss(*args, **kw)
    for kw, text in ((dict(temperature=0.0), "temperature"), (dict(alpha=1.5, labels=lab), "alpha")):
        with pytest.raises(RuntimeError, match=text):
            core.distill_loss(z, ids, top, **kw)
    with pytest.raises(RuntimeError, match="1024"):
        core.distill_loss(z, ids.repeat(1, 300), top.repeat(1, 300))


def test_widths_past_32_bits_are_refused():
    """A vocabulary or a number of entries that 32 bits would cut to a small one is refused, not taken as that."""
    wide = torch.zeros(1, 1, device="cuda").expand(2, 2 ** 32 + 1)
    ids = torch.zeros(1, 1, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="limits"):
        core.distill_loss(wide, ids.expand(2, 3), torch.zeros(2, 3, device="cuda"))
    with pytest.raises(ValueError, match="limits"):
        core.distill_loss(torch.zeros(2, 9, device="cuda"), ids.expand(2, 2 ** 32 + 1), wide)


@pytest.mark.parametrize("go", [1.0, 0.3])
def test_captured_training_step_replays(go):
    z, ids, top, lab = (t.cuda() for t in make(70, 4099, 9, torch.bfloat16, 17))
    outer = torch.tensor(go, device="cuda")

    def step():
        zz = z.detach().requires_grad_(True)
        loss = core.distill_loss(zz, ids, top, labels=lab, alpha=0.4, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss, zz, outer)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dz = step()
    for r in range(4):
        for old, new in zip((z, ids, top, lab), make(70, 4099, 9, torch.bfloat16, 100 + r)):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        wl, wd = step()
        assert torch.equal(loss, wl) and torch.equal(dz, wd), r


def test_two_streams_at_once():
    work = [tuple(t.cuda() for t in make(200, 5000, 8, torch.float32, 20 + s)) for s in range(2)]
    want = [core.distill_loss(z, i, t, labels=y, alpha=0.5) for z, i, t, y in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [None, None]
    for _ in range(3):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                z, i, t, y = work[s]
                got[s] = core.distill_loss(z, i, t, labels=y, alpha=0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("amp", [False, True])
def test_model_distils(amp):
    """OneSdmLM.distill_loss: the loss of its own logits, and a training step whose gradients are those of the same loss put
    together from torch's ops on the same logits."""
    torch.manual_seed(0)
    m = OneSdmLM(211, d=64, layers=2, mlp_f=64, heads=4, n_sub=8, d_a=16, k=4, emb_scale=8.0).cuda()
    g = torch.Generator().manual_seed(3)
    idx = torch.randint(0, 211, (2, 50), generator=g).cuda()
    _, ids, top, lab = (t.cuda() for t in make(100, 211, 7, torch.float32, 21))
    ids, top, lab = ids.view(2, 50, 7), top.view(2, 50, 7), lab.view(2, 50)
    with torch.autocast("cuda", torch.bfloat16, enabled=amp):
        loss = m.distill_loss(idx, ids, top, lab, temperature=2.0, alpha=0.5)
        logits = m(idx)
    assert logits.dtype == (torch.bfloat16 if amp else torch.float32)
    loss.backward()
    rows, grad, lb, _, target, n = reference(logits.detach().cpu().view(100, 211), ids.cpu().view(100, 7), top.cpu().view(100, 7),
                                            lab.cpu().view(100), 2.0, 0.5)
    assert abs(float(loss) - float(rows.sum()) / n) <= float(lb.sum()) / n
    got = {n_: p.grad.clone() for n_, p in m.named_parameters() if p.grad is not None}
    m.zero_grad()
    logits.backward(grad.view(2, 50, 211).to(logits))
    # the two gradients of the logits differ by a rounding of each value: one half step of its type against the other
    rel = 4 * torch.finfo(logits.dtype).eps if amp else 1e-4
    for n_, p in m.named_parameters():
        if p.grad is not None:
            assert float((p.grad - got[n_]).norm()) <= rel * float(p.grad.norm()) + 1e-12, n_


def test_rows_past_32_bits_of_offset():
    """Logits of more than 2^31 elements: the last rows' gradient lies past 32 bits of offset."""
    V, N = 262144, 8200
    z = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    z[-3:] = torch.randn(3, V, generator=torch.Generator().manual_seed(1)).bfloat16().cuda() * 2
    ids = torch.full((N, 2), -1, device="cuda")
    ids[-3:] = torch.tensor([[5, 7], [V - 1, 0], [100, 100]], device="cuda")
    top = torch.tensor([1.0, 2.0], device="cuda").expand(N, 2)
    zz = z.requires_grad_(True)
    loss = core.distill_loss(zz, ids, top)
    dz, = torch.autograd.grad(loss, zz)
    assert not dz[:8].any() and not dz[-20:-3].any()
    rows, grad, lb, gb, _, n = reference(z.detach()[-3:].cpu(), ids[-3:].cpu(), top[-3:].cpu(), None, 1.0, 1.0)
    assert n == 3 and abs(float(loss) - float(rows.sum()) / 3) <= float(lb.sum()) / 3
    err = (dz[-3:].double().cpu() - grad).abs()
    assert bool((err <= gb * 1.01 + 2.0 ** -8 * grad.abs() + 2.0 ** -126).all())
